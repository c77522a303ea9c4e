"""token_log_probs and embed_tokens against plain 64-bit computations.

Tolerances.  A rounding to bf16 is off by at most 2^-8 relative, to fp32 by 2^-24.
Sums of one row: each term e^(x - m) is off by at most 2^-20 relative where it
matters (the argument's rounding, |x - m| < 16, and the exponential's 2^-22), a
thread adds at most 256 terms in order and the tree 12 more, so log s and t / s are
off by at most (256 + 12) 2^-24 + 2^-20 < 2^-15.9 relative to their terms."""

import math

import pytest
import torch

from cyclic_flow_attention import _lib
from cyclic_flow_attention.ops import embed_tokens, token_log_probs

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SUM = 2.0 ** -15.9
BF, F = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _plain(x, tokens, top, ignore=-100):
    """logp, entropy, top values and indices of x (any dtype) in 64 bits."""
    x = x.detach().double()
    m = x.amax(-1, keepdim=True)
    empty = m == -math.inf
    d = torch.where(empty, torch.full_like(x, -math.inf), x - torch.where(empty, 0.0, m))
    s = d.exp().sum(-1, keepdim=True)
    lp = torch.where(empty, d, d - s.log())
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    H = torch.where(x.isnan().any(-1), math.nan, H)
    live = tokens != ignore
    logp = torch.where(live, lp.gather(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None])[..., 0], 0.0)
    order = x.sort(dim=-1, descending=True, stable=True).indices[..., :top]
    return logp, H, lp.gather(-1, order), order, lp, p


def _check(x, tokens, top, grad=True, ignore=-100, seed=0):
    x = x.detach().requires_grad_(grad)
    r = token_log_probs(x, tokens, top=top, ignore_index=ignore)
    logp, H, top_lp, order, lp, p = _plain(x, tokens, top, ignore)
    tol = lambda ref: SUM * (1 + ref.abs().nan_to_num(0, 0, 0)) + 2.0 ** -23 * ref.abs().nan_to_num(0, 0, 0)

    def close(a, b, what):
        same = (a.double() == b) | (a.isnan() & b.isnan())
        bad = ~(same | ((a.double() - b).abs() <= tol(b)))
        assert not bad.any(), (what, a[bad][:5], b[bad][:5])

    close(r.logp, logp, "logp")
    # t / s is a weighted mean of x - m, as large as the entropy or log V
    close(r.entropy, H, "entropy")
    if top:
        assert torch.equal(r.top_tokens, order)
        close(r.top_logp, top_lp, "top_logp")
    else:
        assert r.top_logp is None and r.top_tokens is None
    if grad and tokens.numel():
        g = torch.randn(tokens.shape, generator=_gen(seed + 1), device="cuda")
        h = torch.randn(tokens.shape, generator=_gen(seed + 2), device="cuda")
        dx, = torch.autograd.grad((r.logp, r.entropy), x, (g, h))
        gd = torch.where(tokens != ignore, g, torch.zeros_like(g)).double()[..., None]
        hd = h.double()[..., None]
        inner = torch.where(p > 0, lp, torch.zeros_like(lp)) + H[..., None]
        hit = torch.zeros_like(p).scatter_(-1, tokens.clamp(0, x.shape[-1] - 1)[..., None], 1.0)
        empty = (x.detach().double().amax(-1, keepdim=True) == -math.inf)
        ref = gd * hit - p * (gd + hd * inner)
        ref = torch.where(empty, gd * hit, ref)
        scale = p * (gd.abs() + hd.abs() * (inner.abs() + H[..., None].abs() + 1)) + gd.abs() * hit
        bound = HALF[x.dtype] * 1.01 * ref.abs() + 3 * SUM * scale + 1e-37
        assert dx.dtype == x.dtype and dx.shape == x.shape
        bad = ~((dx.double() - ref).abs() <= bound) & ~(dx.isnan() & ref.isnan())
        assert not bad.any(), (dx[bad][:5], ref[bad][:5])
    return r


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("rows, V, top", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (1, 33, 32), (5, 127, 20),
                                          (2, 640, 32), (257, 1000, 0), (1, 32000, 5), (40, 32003, 20),
                                          (300, 4099, 8), (2, 131072, 32), (1, 262145, 4)])
def test_log_probs_sizes(dtype, rows, V, top):
    x = (torch.randn(rows, V, generator=_gen(V), device="cuda") * 3).to(dtype)
    tokens = torch.randint(V, (rows,), generator=_gen(rows), device="cuda")
    if rows > 2:
        tokens[1] = -100
    _check(x, tokens, top)


@pytest.mark.parametrize("dtype", [BF, F])
def test_log_probs_strides(dtype):
    """Sliced, padded, transposed and expanded logits; rows at every alignment."""
    B, T, V = 3, 5, 515
    big = (torch.randn(B, T + 1, V + 13, generator=_gen(1), device="cuda") * 2).to(dtype)
    tokens = torch.randint(V, (B, T), generator=_gen(2), device="cuda")
    for x in (big[:, :-1, :V], big[:, 1:, 5:V + 5], big[:, 1:, 13:], big[:, ::2, :V][:, :3],
              big.transpose(0, 1)[:T, :, 3:V + 3], big[:1, :T, :V].expand(B, T, V)):
        t = tokens if x.shape[:2] == (B, T) else torch.randint(V, x.shape[:2], generator=_gen(3),
                                                               device="cuda")
        _check(x, t, 4)
    cols = (torch.randn(V, 6, generator=_gen(4), device="cuda")).to(dtype).t()  # last dim strided
    _check(cols, tokens.reshape(-1)[:6], 4)
    x1 = big[0, 0, :V]  # no leading dimension
    _check(x1, tokens[0, 0], 3)
    x4 = big[:, :4, :V].reshape(3, 2, 2, V)
    _check(x4, tokens[:, :4].reshape(3, 2, 2), 3)


def test_log_probs_int32_tokens_and_empty():
    x = torch.randn(4, 100, generator=_gen(0), device="cuda")
    t = torch.randint(100, (4,), generator=_gen(1), device="cuda")
    a, b = token_log_probs(x, t, top=2), token_log_probs(x, t.int(), top=2)
    assert torch.equal(a.logp, b.logp) and torch.equal(a.top_tokens, b.top_tokens)
    e = x[:0].requires_grad_()
    r = token_log_probs(e, t[:0], top=2)
    assert r.logp.shape == (0,) and r.top_tokens.shape == (0, 2)
    g, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), e)
    assert g.shape == (0, 100)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [90, 5000, 40000])
def test_log_probs_masks(dtype, V):
    """-inf masks (also all of a row, all but one), the type's lowest value, NaN,
    +inf, and the token itself masked."""
    x = (torch.randn(9, V, generator=_gen(V), device="cuda") * 3).to(dtype)
    tokens = torch.randint(V, (9,), generator=_gen(1), device="cuda")
    x[1] = -math.inf
    x[2] = -math.inf
    x[2, V - 1] = 1.5
    tokens[2] = V - 1
    x[3, ::2] = -math.inf
    x[4] = torch.finfo(dtype).min
    x[5, 5:] = torch.finfo(dtype).min
    x[6, 3] = math.nan
    x[7, :] = -math.inf
    x[7, 4:V:V // 3] = 0.25
    x[8, 7] = -math.inf
    tokens[8] = 7
    _check(x, tokens, 5)
    top = token_log_probs(x, tokens, top=5)
    assert top.top_tokens[6, 0] == 3 and top.logp[6].isnan() and top.top_logp[6].isnan().all()
    assert torch.equal(top.top_tokens[1].cpu(), torch.arange(5))
    x[6, 3] = math.inf
    r = token_log_probs(x, tokens, top=2)
    assert r.logp[6].isnan() and r.entropy[6].isnan() and r.top_tokens[6, 0] == 3
    assert r.logp[1] == -math.inf and r.entropy[1] == 0 and r.logp[8] == -math.inf
    assert r.entropy[2] == 0 and r.logp[2] == 0


@pytest.mark.parametrize("V", [513, 8192, 70000])
def test_log_probs_ties_and_runs(V):
    """Equal values, both zeros, sorted rows and all large values side by side:
    the order is by value, then lowest index."""
    x = torch.zeros(6, V, device="cuda")
    x[1] = torch.where(torch.arange(V, device="cuda") % 2 == 0, -0.0, 0.0)
    x[2] = torch.arange(V, device="cuda") / V
    x[3] = -torch.arange(V, device="cuda") / V
    at = torch.arange(V, device="cuda")
    x[4] = ((at // 8) % 512 < 5).float() + torch.rand(V, generator=_gen(3), device="cuda") * 0.5
    x[5] = torch.randint(3, (V,), generator=_gen(4), device="cuda").float()
    tokens = torch.randint(V, (6,), generator=_gen(5), device="cuda")
    for dtype in (F, BF):
        for top in (1, 20, 32):
            _check(x.to(dtype), tokens, top)


def test_log_probs_bad_token_is_reported():
    _lib.device_error()
    x = torch.randn(3, 50, generator=_gen(0), device="cuda").requires_grad_()
    r = token_log_probs(x, torch.tensor([4, 50, -3], device="cuda"))
    assert r.logp[0].isfinite() and r.logp[1:].isnan().all() and r.entropy.isfinite().all()
    g, = torch.autograd.grad(r.logp, x, torch.ones(3, device="cuda"))
    assert (g[1:] == 0).all() and (g[0] != 0).any()
    assert _lib.device_error() == 3 and _lib.device_error() == 0


def test_log_probs_one_gradient_at_a_time_and_twice():
    x = torch.randn(7, 333, generator=_gen(0), device="cuda").requires_grad_()
    t = torch.randint(333, (7,), generator=_gen(1), device="cuda")
    r = token_log_probs(x, t, top=3)
    assert not r.top_logp.requires_grad
    a, = torch.autograd.grad(r.logp.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(r.entropy.sum(), x, retain_graph=True)
    c, = torch.autograd.grad(r.logp.sum() + r.entropy.sum(), x)
    torch.testing.assert_close(a + b, c, rtol=1e-5, atol=1e-6)
    y = x.detach().double().cpu().requires_grad_()
    lp = torch.log_softmax(y, -1)
    ref, = torch.autograd.grad(lp.gather(-1, t.cpu()[:, None]).sum(), y)
    assert (a.double().cpu() - ref).abs().max() < 2.0 ** -14


def test_log_probs_gradient_by_differences():
    """(f(x + e) - f(x - e)) / 2e of the 64-bit formula against the kernel's gradient."""
    x = torch.randn(2, 20, generator=_gen(0), device="cuda")
    t = torch.randint(20, (2,), generator=_gen(1), device="cuda")
    xr = x.clone().requires_grad_()
    r = token_log_probs(xr, t)
    g, = torch.autograd.grad((r.logp * 0.7 + r.entropy * 1.3).sum(), xr)
    e = 1e-5
    for i in range(2):
        for j in range(20):
            d = torch.zeros(2, 20, dtype=torch.float64, device="cuda")
            d[i, j] = e
            f = [(_plain(x.double() + s * d, t, 1)[0] * 0.7 + _plain(x.double() + s * d, t, 1)[1] * 1.3).sum()
                 for s in (1, -1)]
            assert abs(float(f[0] - f[1]) / (2 * e) - float(g[i, j])) < 1e-4


def test_log_probs_offsets_past_32_bits():
    """Rows whose first element lies beyond 2^32 elements."""
    stride = 2_300_000_008
    buf = torch.empty(2 * stride + 4096, device="cuda", dtype=BF)
    x = buf.as_strided((3, 1000), (stride, 1))
    x.copy_((torch.randn(3, 1000, generator=_gen(0), device="cuda")).to(BF))
    t = torch.randint(1000, (3,), generator=_gen(1), device="cuda")
    a, b = token_log_probs(x, t, top=4), token_log_probs(x.clone(), t, top=4)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_log_probs_stream_graph_and_repeat():
    """Another stream, a captured and replayed call with new inputs, and the same
    bits twice."""
    x = torch.randn(64, 8000, generator=_gen(0), device="cuda").to(BF).requires_grad_()
    t = torch.randint(8000, (64,), generator=_gen(1), device="cuda")
    g = torch.randn(64, generator=_gen(2), device="cuda")

    def step():
        r = token_log_probs(x, t, top=6)
        dx, = torch.autograd.grad((r.logp, r.entropy), x, (g, g))
        # (results that keep their autograd graph alive would tie the leaf to this stream)
        return [v.detach() for v in r] + [dx]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn(64, 8000, generator=_gen(3), device="cuda"))
    t.copy_(torch.randint(8000, (64,), generator=_gen(4), device="cuda"))
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


# ------------------------------------------------------------------- embedding
def _embed_check(tokens, weight, scale=1.0, padding_idx=None, seed=0):
    w = weight.detach().requires_grad_()
    out = embed_tokens(tokens, w, scale=scale, padding_idx=padding_idx)
    ref = w.detach()[tokens.long()].double() * scale
    half = HALF[w.dtype] * 1.01
    assert out.dtype == w.dtype
    assert ((out.double() - ref).abs() <= half * ref.abs() + 2.0 ** -23 * ref.abs()).all()
    dout = torch.randn(out.shape, generator=_gen(seed), device="cuda").to(w.dtype)
    dw, = torch.autograd.grad(out, w, dout)
    flat, d = tokens.long().reshape(-1), dout.reshape(-1, w.shape[1]).double()
    sums = torch.zeros(w.shape, dtype=torch.float64, device="cuda").index_add_(0, flat, d) * scale
    mags = torch.zeros(w.shape, dtype=torch.float64, device="cuda").index_add_(0, flat, d.abs())
    if padding_idx is not None:
        sums[padding_idx] = 0
        mags[padding_idx] = 0
    count = torch.bincount(flat, minlength=w.shape[0]).double()[:, None]
    bound = half * sums.abs() + (count + 2) * 2.0 ** -24 * mags * abs(scale)
    bad = ~((dw.double() - sums).abs() <= bound)
    assert not bad.any(), (bad.nonzero()[:5], dw[bad][:5], sums[bad][:5])
    dw2, = torch.autograd.grad(embed_tokens(tokens, w, scale=scale, padding_idx=padding_idx), w, dout)
    assert torch.equal(dw, dw2)


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("N, V, D", [(1, 1, 1), (1, 300, 8), (31, 2, 3), (32, 5, 16), (33, 7, 129),
                                     (1000, 255, 64), (1000, 256, 63), (4097, 257, 40), (5000, 70000, 24),
                                     (9000, 3, 520), (2048, 32000, 1024), (700, 16777300, 4)])
def test_embedding_sizes(dtype, N, V, D):
    w = torch.randn(V, D, generator=_gen(V), device="cuda").to(dtype)
    tokens = torch.randint(V, (N,), generator=_gen(N), device="cuda")
    _embed_check(tokens, w, scale=0.5 if N % 2 else 1.7)


@pytest.mark.parametrize("dtype", [BF, F])
def test_embedding_runs(dtype):
    """One id for all tokens, runs that end at, before and after the pieces' ends,
    first and last ids, padding rows, shapes and int32."""
    V, D = 50, 72
    w = torch.randn(V, D, generator=_gen(0), device="cuda").to(dtype)
    _embed_check(torch.full((100000,), 7, device="cuda"), w)
    for run in (1, 31, 32, 33, 63, 64, 65, 96, 1000):
        _embed_check(torch.arange(40 * run, device="cuda") // run % V, w, seed=run)
    t = torch.randint(V, (6, 7, 11), generator=_gen(1), device="cuda")
    t[0] = 0
    t[1] = V - 1
    _embed_check(t, w, padding_idx=0)
    _embed_check(t.int(), w, padding_idx=-1)
    _embed_check(t.transpose(0, 2), w)
    _embed_check(torch.full((3000,), 4, device="cuda"), w, padding_idx=4)


@pytest.mark.parametrize("N, V", [(131072, 90000), (131073, 90000), (200003, 300), (300000, 16777300)])
def test_embedding_many_tokens(N, V):
    """Both sides of the number of tokens that one cluster sorts, with runs, a
    padding row and tokens outside the vocabulary."""
    w = torch.randn(V, 4, generator=_gen(0), device="cuda")
    t = torch.randint(V, (N,), generator=_gen(1), device="cuda")
    t[N // 3: N // 2] = V - 1
    t[::7] = 5
    _embed_check(t, w, padding_idx=5)
    w = w.requires_grad_()
    bad = t.clone()
    bad[::5], bad[1::11] = -1, V
    d = torch.randn(N, 4, generator=_gen(2), device="cuda")
    _lib.device_error()
    g, = torch.autograd.grad(embed_tokens(bad, w), w, d)
    ok = (bad >= 0) & (bad < V)
    want, = torch.autograd.grad(embed_tokens(bad[ok], w), w, d[ok])
    assert torch.equal(g, want)  # the dropped entries come last: the same sums
    assert _lib.device_error() == 3


def test_embedding_misaligned_and_strided_table():
    big = torch.randn(40, 70, generator=_gen(0), device="cuda")
    t = torch.randint(40, (500,), generator=_gen(1), device="cuda")
    for w in (big[:, 1:65], big.t()[:40, :40], torch.randn(40 * 64 + 1, device="cuda")[1:].view(40, 64)):
        _embed_check(t % w.shape[0], w)
        _embed_check(t % w.shape[0], w.to(BF))


def test_embedding_empty_bad_tokens_and_gradient_strides():
    w = torch.randn(20, 8, generator=_gen(0), device="cuda").requires_grad_()
    out = embed_tokens(torch.zeros(0, 3, dtype=torch.long, device="cuda"), w)
    assert out.shape == (0, 3, 8)
    g, = torch.autograd.grad(out.sum(), w)
    assert (g == 0).all() and g.shape == w.shape
    _lib.device_error()
    t = torch.tensor([3, 20, -1, 5, -100, 3], device="cuda")
    out = embed_tokens(t, w)
    assert (out[[1, 2, 4]] == 0).all() and torch.equal(out[3], w[5])
    dout = torch.randn(8, 6, generator=_gen(1), device="cuda").t()  # a strided gradient
    g, = torch.autograd.grad(out, w, dout)
    ref = torch.zeros(20, 8, device="cuda")
    ref[3], ref[5] = dout[0] + dout[5], dout[3]
    assert torch.equal(g, ref)
    assert _lib.device_error() == 3


def test_embedding_offsets_past_32_bits():
    """A table of more than 2^32 elements, forward and gradient."""
    V, D = 2_200_000, 2048
    w = torch.zeros(V, D, device="cuda", dtype=BF)
    t = torch.tensor([V - 1, 5, V - 2, V - 1, 2_097_153], device="cuda")
    w[t] = torch.randn(5, D, generator=_gen(0), device="cuda").to(BF)
    w.requires_grad_()
    out = embed_tokens(t, w)
    assert torch.equal(out, w.detach()[t])
    dout = torch.randn(5, D, generator=_gen(1), device="cuda").to(BF)
    g, = torch.autograd.grad(out, w, dout)
    assert torch.equal(g[V - 2], dout[2]) and torch.equal(g[5], dout[1])
    assert torch.equal(g[V - 1], (dout[0].float() + dout[3].float()).to(BF))
    assert torch.equal(g[2_097_153], dout[4])
    assert int(torch.count_nonzero(g)) == int(torch.count_nonzero(g[t[1:]]))


def test_embedding_stream_and_graph():
    w = torch.randn(3000, 64, generator=_gen(0), device="cuda").requires_grad_()
    t = torch.randint(3000, (5000,), generator=_gen(1), device="cuda")
    d = torch.randn(5000, 64, generator=_gen(2), device="cuda")
    step = lambda: [(o := embed_tokens(t, w, 2.0, 3)).detach(), torch.autograd.grad(o, w, d)[0]]
    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    t.copy_(torch.randint(40, (5000,), generator=_gen(3), device="cuda"))
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))

"""residual_norm against plain 64-bit computations.

Tolerances.  Rounding: bf16 2^-8, fp32 2^-24 relative.  Sums of squares and dot
products of a row: 8 terms in order per thread and a tree of at most 10, each
2^-24, and the sigmoid's and reciprocal root's few ulp: 2^-18 relative to the terms
covers them.  Column sums: at most 2000 rows in order, 2000 2^-24 < 2^-13 of the
sum of magnitudes."""

import pytest
import torch

from cyclic_flow_attention.ops import residual_norm

pytestmark = pytest.mark.gpu
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
ROW, COL = 2.0 ** -18, 2.0 ** -13
BF, F = torch.bfloat16, torch.float32
EPS = 1e-6


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(shape, dtype, post, gate, scale, seed=0, wdtype=F):
    g = _gen(seed)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    D = shape[-1]
    return dict(
        x=(2 * n(*shape)).to(dtype), y=n(*shape).to(dtype), weight=(1 + 0.3 * n(D)).to(wdtype),
        post_weight=(1 + 0.3 * n(D)).to(wdtype) if post else None,
        gate=n(*shape).to(dtype) if gate else None,
        scale={"none": None, "number": -0.7, "vector": (0.5 + n(D)).to(wdtype)}[scale])


def _check(ins, grad=True, dx_given=True, dh_given=True, seed=1):
    dtype = ins["x"].dtype
    half, D = HALF[dtype] * 1.01, ins["x"].shape[-1]
    leaf = {k: (t.detach().requires_grad_(grad) if isinstance(t, torch.Tensor) else t)
            for k, t in ins.items()}
    xn, h = residual_norm(leaf["x"], leaf["y"], leaf["weight"], leaf["post_weight"], leaf["gate"],
                          leaf["scale"], EPS)
    assert xn.dtype == h.dtype == dtype and xn.shape == h.shape == ins["x"].shape
    q = {k: (t.detach().double() if isinstance(t, torch.Tensor) else t) for k, t in ins.items()}
    y, post = q["y"], q["post_weight"]
    ny = (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() if post is not None else 1.0
    yh = y / ny
    z = yh * post if post is not None else yh
    sg = torch.sigmoid(q["gate"]) if q["gate"] is not None else torch.ones_like(y)
    sc = 1.0 if q["scale"] is None else q["scale"]
    u = sc * sg * z
    ref = q["x"] + u
    err = (xn.double() - ref).abs()
    assert (err <= half * ref.abs() + ROW * (q["x"].abs() + u.abs())).all()
    # the norm acts on the stream as the kernel rounded it
    t = xn.detach().double()
    nt = (t.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    th = t / nt
    ref = th * q["weight"]
    assert ((h.double() - ref).abs() <= (half + ROW) * ref.abs()).all()
    if not grad:
        return xn, h
    dxn = torch.randn(xn.shape, generator=_gen(seed), device="cuda").to(dtype)
    dh = torch.randn(xn.shape, generator=_gen(seed + 1), device="cuda").to(dtype)
    outs = ([xn] if dx_given else []) + ([h] if dh_given else [])
    gos = ([dxn] if dx_given else []) + ([dh] if dh_given else [])
    names = [k for k, v in leaf.items() if isinstance(v, torch.Tensor) and (dh_given or k != "weight")]
    got = dict(zip(names, torch.autograd.grad(outs, [leaf[k] for k in names], gos)))
    a = dxn.double() if dx_given else torch.zeros_like(t)
    b = dh.double() if dh_given else torch.zeros_like(t)
    bw = b * q["weight"]
    dot = (bw * th).mean(-1, keepdim=True)
    dt = a + (bw - th * dot) / nt
    mt = a.abs() + (bw.abs() + th.abs() * (bw * th).abs().mean(-1, keepdim=True)) / nt
    dz, mz = dt * sc * sg, mt * (sg * abs(sc) if not isinstance(sc, torch.Tensor) else sg * sc.abs())
    dy, my = dz, mz
    if post is not None:
        w = dz * post
        mw = mz * post.abs()
        dy = (w - yh * (w * yh).mean(-1, keepdim=True)) / ny
        my = (mw + yh.abs() * (mw * yh.abs()).mean(-1, keepdim=True)) / ny
    asc = sc.abs() if isinstance(sc, torch.Tensor) else abs(sc)
    rowwise = {"x": (dt, mt), "y": (dy, my),
               "gate": (dt * sc * z * sg * (1 - sg), mt * asc * z.abs() * sg * (1 - sg))}
    flat = lambda v: v.reshape(-1, D)
    column = {"weight": (b * th, b.abs() * th.abs()), "post_weight": (dz * yh, mz * yh.abs()),
              "scale": (dt * sg * z, mt * sg * z.abs())}
    for k, g in got.items():
        assert g.dtype == leaf[k].dtype and g.shape == leaf[k].shape
        if k in rowwise:
            r, m = rowwise[k]
            bound = half * r.abs() + 4 * ROW * m
        else:
            r, m = (flat(v).sum(0) for v in column[k])
            bound = HALF[leaf[k].dtype] * 1.01 * r.abs() + COL * m
        bad = ~((g.double() - r).abs() <= bound)
        assert not bad.any(), (k, g[bad][:5], r[bad][:5])
    return xn, h


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("rows, D", [(1, 1), (3, 2), (5, 7), (2, 8), (33, 100), (17, 256), (9, 257), (300, 1024),
                                     (7, 1531), (40, 2048), (5, 4099), (3, 8191), (4, 8192), (2000, 64)])
def test_sizes(dtype, rows, D):
    _check(_inputs((rows, D), dtype, False, False, "none"))
    _check(_inputs((rows, D), dtype, True, True, "vector"))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("scale", ["none", "number", "vector"])
def test_forms(dtype, post, gate, scale):
    _check(_inputs((2, 21, 136), dtype, post, gate, scale))
    _check(_inputs((2, 21, 136), dtype, post, gate, scale), dx_given=False)
    _check(_inputs((2, 21, 136), dtype, post, gate, scale), dh_given=False)
    _check(_inputs((45, 130), dtype, post, gate, scale, wdtype=BF), grad=False)
    _check(_inputs((45, 130), dtype, post, gate, scale, wdtype=BF))


@pytest.mark.parametrize("dtype", [BF, F])
def test_norm_alone(dtype):
    x = torch.randn(50, 96, generator=_gen(0), device="cuda").to(dtype).requires_grad_()
    w = (1 + torch.randn(96, generator=_gen(1), device="cuda")).requires_grad_()
    xn, h = residual_norm(x, None, w, eps=EPS)
    assert xn is x
    t = x.detach().double()
    n = (t.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    ref = t / n * w.detach().double()
    assert ((h.double() - ref).abs() <= (HALF[dtype] * 1.01 + ROW) * ref.abs()).all()
    dh = torch.randn(h.shape, generator=_gen(2), device="cuda").to(dtype)
    dx, dw = torch.autograd.grad(h, (x, w), dh)
    b = dh.double() * w.detach().double()
    r = (b - t / n * (b * t / n).mean(-1, keepdim=True)) / n
    m = (b.abs() + (t / n).abs() * (b * t / n).abs().mean(-1, keepdim=True)) / n
    assert ((dx.double() - r).abs() <= HALF[dtype] * 1.01 * r.abs() + 4 * ROW * m).all()
    assert ((dw.double() - (dh.double() * t / n).sum(0)).abs() <= COL * (dh.double() * t / n).abs().sum(0)).all()


@pytest.mark.parametrize("dtype", [BF, F])
def test_strides(dtype):
    """Column views of a packed projection, odd offsets, transposed and expanded inputs."""
    B, T, D = 3, 10, 64
    packed = torch.randn(B, T, 5 * D + 3, generator=_gen(0), device="cuda").to(dtype)
    base = _inputs((B, T, D), dtype, True, True, "vector")
    for lo in (0, 1, 8):
        ins = dict(base, y=packed[..., lo:lo + D], gate=packed[..., 2 * D + lo:3 * D + lo])
        _check(ins)
    _check(dict(base, x=packed.transpose(0, 1)[..., :D].reshape(T, B, D).transpose(0, 1)))
    _check(dict(base, gate=packed[:, :1, :D].expand(B, T, D)))
    _check(dict(base, x=torch.randn(D, B, T, generator=_gen(3), device="cuda").to(dtype).permute(1, 2, 0)))


def test_broadcast_gate_gradient():
    """A gate of one row per sequence, expanded by the caller: its gradient sums
    over the tokens."""
    ins = _inputs((2, 9, 40), F, False, False, "none")
    g1 = torch.randn(2, 1, 40, generator=_gen(5), device="cuda").requires_grad_()
    g2 = g1.detach().expand(2, 9, 40).contiguous().requires_grad_()
    out = []
    for g in (g1.expand(2, 9, 40), g2):
        xn, h = residual_norm(ins["x"], ins["y"], ins["weight"], gate=g)
        out.append((xn * 0.3 + h * h).sum())
    a, = torch.autograd.grad(out[0], g1)
    b, = torch.autograd.grad(out[1], g2)
    torch.testing.assert_close(a, b.sum(1, keepdim=True), rtol=1e-5, atol=1e-5)


def test_gradient_by_differences():
    ins = _inputs((2, 6), F, True, True, "vector")
    leaf = {k: t.clone().requires_grad_() for k, t in ins.items()}
    c = torch.randn(2, 2, 6, generator=_gen(9), device="cuda").double()

    def f(v):
        y, post = v["y"], v["post_weight"]
        z = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * post
        xn = v["x"] + v["scale"] * torch.sigmoid(v["gate"]) * z
        h = xn / (xn.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * v["weight"]
        return (c[0] * xn + c[1] * h).sum()

    xn, h = residual_norm(leaf["x"], leaf["y"], leaf["weight"], leaf["post_weight"], leaf["gate"],
                          leaf["scale"], EPS)
    grads = torch.autograd.grad((xn, h), list(leaf.values()), (c[0].float(), c[1].float()))
    base = {k: t.double() for k, t in ins.items()}
    for (k, t), g in zip(leaf.items(), grads):
        for i in range(t.numel()):
            d = torch.zeros(t.numel(), dtype=torch.float64, device="cuda")
            d[i] = 1e-5
            d = d.view(t.shape)
            num = (f(dict(base, **{k: base[k] + d})) - f(dict(base, **{k: base[k] - d}))) / 2e-5
            assert abs(float(num) - float(g.reshape(-1)[i])) < 1e-4 * (1 + abs(float(num))), (k, i)


def test_zero_rows_empty_and_special_values():
    x = torch.zeros(4, 48, device="cuda", requires_grad=True)
    y = torch.zeros(4, 48, device="cuda", requires_grad=True)
    w = torch.ones(48, device="cuda", requires_grad=True)
    xn, h = residual_norm(x, y, w, post_weight=w)
    assert (xn == 0).all() and (h == 0).all()
    g = torch.autograd.grad(h.sum(), (x, y, w))
    assert all(t.isfinite().all() for t in g)
    gate = torch.full((4, 48), -200.0, device="cuda")
    gate[:, ::2] = 200.0
    y = torch.ones(4, 48, device="cuda", requires_grad=True)
    gate.requires_grad_()
    xn, h = residual_norm(x, y, w, gate=gate)
    assert (xn[:, ::2] == 1).all() and (xn[:, 1::2] == 0).all()
    assert all(t.isfinite().all() for t in torch.autograd.grad((xn.sum() + h.sum()), (x, y, gate, w)))
    z = torch.zeros(0, 48, device="cuda", requires_grad=True)
    xn, h = residual_norm(z, torch.zeros(0, 48, device="cuda"), w)
    gz, gw = torch.autograd.grad(h.sum(), (z, w))
    assert gz.shape == (0, 48) and (gw == 0).all()
    x = torch.ones(3, 16, device="cuda")
    x[1, 3] = float("nan")
    _, h = residual_norm(x, None, torch.ones(16, device="cuda"))
    assert h[1].isnan().all() and h[0].isfinite().all() and h[2].isfinite().all()


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("D", [64, 67, 1024])
@pytest.mark.parametrize("post, gate, scale", [(False, False, "none"), (False, True, "number"),
                                               (True, False, "vector"), (True, True, "number")])
def test_infinities_follow_the_formula(dtype, D, post, gate, scale):
    """Infinite and overflowing entries give the formula's infinities, zeros and NaN
    in fp32, and leave the other rows alone.  Tolerance: one step of x's type on x'
    (it may round to the neighbour), and on h, which is the formula of the x' returned:
    where x and z cancel, fp32's 2^-24 |x| is any multiple of x' and so of h."""
    ins = _inputs((7, D), dtype, post, gate, scale)
    inf = float("inf")
    ins["x"][0, 3], ins["x"][1, 5] = inf, -inf
    ins["y"][2, 4], ins["y"][3, 6] = inf, -inf
    ins["y"][4, 1] = 3e38
    if gate:
        ins["gate"][5, 2], ins["gate"][5, 7], ins["gate"][2, 9] = inf, -inf, -inf
    xn, h = residual_norm(ins["x"], ins["y"], ins["weight"], ins["post_weight"], ins["gate"],
                          ins["scale"], EPS)
    z = ins["y"].float()
    if post:
        z = z * torch.rsqrt(z.pow(2).mean(-1, keepdim=True) + EPS) * ins["post_weight"]
    if gate:
        z = z * torch.sigmoid(ins["gate"].float())
    x = (ins["x"].float() + z * (1.0 if ins["scale"] is None else ins["scale"])).to(dtype)
    f = xn.float()
    n = (f * torch.rsqrt(f.pow(2).mean(-1, keepdim=True) + EPS) * ins["weight"]).to(dtype)
    step = 2 * HALF[dtype] if dtype == BF else 2.0 ** -18
    for got, ref, near in ((xn, x, 4), (h, n, 0)):
        assert torch.equal(got.isnan(), ref.isnan())
        keep = ~ref.isnan()
        g, r = got.double()[keep], ref.double()[keep]
        same = g == r
        assert (same | ((g - r).abs() <= 1.01 * step * (r.abs() + near))).all()


def test_offsets_past_32_bits():
    stride = 2_300_000_008
    buf = torch.empty(2 * stride + 4096, device="cuda", dtype=BF)
    x = buf.as_strided((3, 512), (stride, 1))
    x.copy_(torch.randn(3, 512, generator=_gen(0), device="cuda").to(BF))
    w = torch.ones(512, device="cuda")
    a = residual_norm(x, x, w)
    b = residual_norm(x.clone(), x.clone(), w)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_stream_graph_and_repeat():
    ins = _inputs((700, 320), BF, True, True, "vector")
    leaf = {k: t.requires_grad_() for k, t in ins.items()}
    d = torch.randn(700, 320, generator=_gen(2), device="cuda").to(BF)

    def step():
        xn, h = residual_norm(leaf["x"], leaf["y"], leaf["weight"], leaf["post_weight"], leaf["gate"],
                              leaf["scale"])
        return [xn.detach(), h.detach(), *torch.autograd.grad((xn, h), list(leaf.values()), (d, d))]

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
        leaf["x"].copy_(torch.randn(700, 320, generator=_gen(3), device="cuda"))
    graph.replay()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_aliased_inputs():
    """One tensor as stream, branch and gate: its gradient is the sum of the three."""
    x = torch.randn(20, 64, generator=_gen(0), device="cuda").requires_grad_()
    w = torch.ones(64, device="cuda")
    xn, h = residual_norm(x, x, w, gate=x)
    a, = torch.autograd.grad((xn * 0.5 + h).sum(), x)
    xs = [x.detach().clone().requires_grad_() for _ in range(3)]
    xn, h = residual_norm(xs[0], xs[1], w, gate=xs[2])
    b = sum(torch.autograd.grad((xn * 0.5 + h).sum(), xs))
    torch.testing.assert_close(a, b, rtol=1e-5, atol=1e-6)
    xn, h = residual_norm(x, x, w)
    c, = torch.autograd.grad(xn.sum(), x)
    assert torch.equal(c, torch.full_like(c, 2.0))


@pytest.mark.parametrize("width", [1024, 514, 77])
@pytest.mark.parametrize("gate", [False, True])
def test_bf16_stream_is_the_exact_sums_rounding(width, gate):
    """x' in bf16 equals the 64-bit sum rounded to fp32 and then to bf16.  The branch is
    exact to 2^-38 without a gate and 2^-28 with one, relative to |x'| at worst 2^4
    times more; an entry moves when that straddles a rounding border of spacing 2^-8:
    at most 2^-26 and 2^-16 of the 2^18 entries, 0 and a few."""
    ins = _inputs((2 ** 18 // width, width), BF, True, gate, "vector", seed=7)
    xn, _ = residual_norm(ins["x"], ins["y"], ins["weight"], ins["post_weight"], ins["gate"],
                          ins["scale"], EPS)
    y = ins["y"].double()
    u = y / (y.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * ins["post_weight"].double()
    u = u * ins["scale"].double()
    if gate:
        u = u * torch.sigmoid(ins["gate"].double())
    ref = (ins["x"].double() + u).float().to(BF)
    assert int((xn != ref).sum()) <= (4 if gate else 0)

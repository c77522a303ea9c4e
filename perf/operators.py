"""Timed passes of the language-model operators around the CyFA layer.

Four operators, each with its plain form in elementary torch operations and its
definition in 64 bits:

* ``logprobs``  token log probabilities with entropy and top alternatives
* ``embed``     scaled embedding lookup, gradient summed in token order
* ``norm``      residual add with gate, scale and the norms before and after it
* ``newton``    Newton-Schulz orthogonalisation of a matrix update

``run`` takes the plain form while ``own`` is false and the package's operators
while it is true.
"""

import math
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
# quintic Newton-Schulz: X <- a X + (b A + c A A) X with A = X X^T
_QUINTIC = (3.4445, -4.7750, 2.0315)
_STEPS = 5
_NS_EPS = 1e-7
_NORM_EPS = 1e-6
_IGNORE = -100


# ----------------------------------------------------------------- the cases
def listed():
    lp = dict(op="logprobs", strided=False, masked=False)
    em = dict(op="embed", padding=False)
    nm = dict(op="norm")
    ns = dict(op="newton")
    return [
        # one sequence being decoded, its alternatives shown to the user: latency
        lp | dict(name="logprobs_decode_1", batch=1, tokens=1, vocab=32000, dtype="bf16", top=5,
                  grad=False),
        # a decode step of the whole serving batch under a vocabulary mask
        lp | dict(name="logprobs_decode_256", batch=256, tokens=1, vocab=32000, dtype="bf16",
                  top=20, grad=False, masked=True),
        # the loss of a training step (8 sequences of 2048 tokens) and its gradient
        lp | dict(name="logprobs_train", batch=8, tokens=2048, vocab=32000, dtype="bf16", top=0,
                  grad=True),
        # fp32 logits of all positions but the last, odd vocabulary: a policy update
        lp | dict(name="logprobs_odd_f32", batch=8, tokens=129, vocab=50021, dtype="f32", top=3,
                  grad=True, strided=True),
        # one decode step's lookup: latency
        em | dict(name="embed_decode_256", count=256, vocab=32000, width=1024, dtype="bf16",
                  grad=False),
        # the lookup of a training step and the gradient of the whole table
        em | dict(name="embed_train", count=16384, vocab=32000, width=1024, dtype="bf16",
                  grad=True),
        # a large fp32 table of odd width, a tenth of the tokens padding
        em | dict(name="embed_odd_f32", count=30011, vocab=100003, width=1001, dtype="f32",
                  grad=True, padding=True),
        # residual add and norm of one decode step: latency
        nm | dict(name="norm_decode_256", rows=256, width=1024, dtype="bf16", post=False,
                  gate=False, scale="none", grad=False),
        # a block's residual add and norm in a training step, with gradients
        nm | dict(name="norm_train", rows=16384, width=1024, dtype="bf16", post=False, gate=False,
                  scale="none", grad=True),
        # norms on both sides, gate and per-channel scale, odd fp32 sizes
        nm | dict(name="norm_sandwich_odd_f32", rows=4099, width=1531, dtype="f32", post=True,
                  gate=True, scale="vector", grad=True),
        # a few small fp32 matrices of odd shape: launches and latency
        ns | dict(name="newton_small_odd", count=4, m=127, n=509, dtype="f32"),
        # the MLP matrices of 24 layers, as an optimiser's step takes them
        ns | dict(name="newton_mlp", count=24, m=2816, n=1024, dtype="bf16"),
    ]


def _spread(rng, low, high):
    """A whole number, spread evenly over the logarithm of [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["logprobs", "embed", "norm", "newton"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "logprobs":
        vocab = _spread(rng, 128, 131072)
        top = rng.choice([0, 1, 5, 20])
        grad = rng.random() < 0.5
        # a sorted row of the plain form costs far more than a summed one
        limit = (1 << 25) if top else (1 << 28)
        rows = _spread(rng, 1, max(1, min(16384, limit // vocab)))
        batch = rng.choice([b for b in (1, 2, 4, 8) if b <= rows])
        return dict(op=op, batch=batch, tokens=max(1, rows // batch), vocab=vocab, dtype=dtype,
                    top=min(top, vocab), grad=grad, strided=rng.random() < 0.4,
                    masked=rng.random() < 0.3)
    if op == "embed":
        return dict(op=op, count=_spread(rng, 1, 32768), vocab=_spread(rng, 128, 65536),
                    width=_spread(rng, 64, 2048), dtype=dtype, grad=rng.random() < 0.7,
                    padding=rng.random() < 0.4)
    if op == "norm":
        return dict(op=op, rows=_spread(rng, 1, 16384), width=_spread(rng, 32, 4096), dtype=dtype,
                    post=rng.random() < 0.5, gate=rng.random() < 0.5,
                    scale=rng.choice(["none", "number", "vector"]), grad=rng.random() < 0.7)
    return dict(op=op, count=_spread(rng, 1, 16), m=_spread(rng, 16, 2048), n=_spread(rng, 16, 2048),
                dtype=dtype)


# ----------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    s = {"case": case}
    if case["op"] == "logprobs":
        B, T, V = case["batch"], case["tokens"], case["vocab"]
        base = (normal(B, T + 1 if case["strided"] else T, V) * 2.5).to(dt)
        x = base[:, :T]
        tokens = (uniform(B, T) * V).long().clamp_(max=V - 1)
        if case["masked"]:
            kept = x.gather(2, tokens[..., None])
            x.masked_fill_(uniform(V) < 0.3, -math.inf)
            x.scatter_(2, tokens[..., None], kept)
        if case["grad"]:
            # a tenth of the positions carry no loss
            tokens.masked_fill_(uniform(B, T) < 0.1, _IGNORE)
            s["d_logp"] = normal(B, T)
            s["d_entropy"] = normal(B, T) * 0.1
        s["logits"] = x.detach().requires_grad_(case["grad"])
        s["tokens"] = tokens
    elif case["op"] == "embed":
        N, V, D = case["count"], case["vocab"], case["width"]
        # ranks fall off as 1/r, as words do; the order of the ids is shuffled
        rank = torch.exp(uniform(N) * math.log(V)).long().clamp_(1, V) - 1
        tokens = torch.randperm(V, generator=gen, device="cuda")[rank]
        if case["padding"]:
            tokens.masked_fill_(uniform(N) < 0.1, 0)
        s["tokens"] = tokens
        s["weight"] = (normal(V, D) * 0.02).to(dt).requires_grad_(case["grad"])
        s["scale"] = math.sqrt(D)
        if case["grad"]:
            s["d_out"] = normal(N, D).to(dt)
    elif case["op"] == "norm":
        N, D, grad = case["rows"], case["width"], case["grad"]
        s["x"] = (normal(N, D) * 2).to(dt).requires_grad_(grad)
        s["y"] = normal(N, D).to(dt).requires_grad_(grad)
        s["weight"] = (1 + 0.1 * normal(D)).requires_grad_(grad)
        s["post"] = (1 + 0.1 * normal(D)).requires_grad_(grad) if case["post"] else None
        s["gate"] = normal(N, D).to(dt).requires_grad_(grad) if case["gate"] else None
        s["scale"] = {"none": None, "number": 0.5,
                      "vector": (0.5 + 0.1 * normal(D)).requires_grad_(grad)}[case["scale"]]
        if grad:
            s["d_x"] = normal(N, D).to(dt)
            s["d_h"] = normal(N, D).to(dt)
    else:
        L, m, n = case["count"], case["m"], case["n"]
        # a gradient: a few strong directions over noise
        r = max(1, min(m, n) // 16)
        g = normal(L, m, r) @ (normal(L, r, n) * 0.2) + normal(L, m, n) * 0.1
        s["g"] = (g * 1e-3).to(dt)
    return s


# ----------------------------------------------------------------- the passes
def _package():
    root = os.path.join(os.getcwd(), "cyfa-jittor_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cyclic_flow_attention import ops
    return ops


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    ops, case = _package(), s["case"]
    if case["op"] == "logprobs":
        r = ops.token_log_probs(s["logits"], s["tokens"], top=case["top"], ignore_index=_IGNORE)
        out = {"logp": r.logp, "entropy": r.entropy}
        if case["top"]:
            out |= {"top_logp": r.top_logp, "top_tokens": r.top_tokens}
        if case["grad"]:
            out["d_logits"], = torch.autograd.grad(
                (r.logp, r.entropy), (s["logits"],), (s["d_logp"], s["d_entropy"]))
        return out
    if case["op"] == "embed":
        h = ops.embed_tokens(s["tokens"], s["weight"], scale=s["scale"],
                             padding_idx=0 if case["padding"] else None)
        out = {"h": h}
        if case["grad"]:
            out["d_weight"], = torch.autograd.grad((h,), (s["weight"],), (s["d_out"],))
        return out
    if case["op"] == "norm":
        x, h = ops.residual_norm(s["x"], s["y"], s["weight"], post_weight=s["post"],
                                 gate=s["gate"], scale=s["scale"], eps=_NORM_EPS)
        out = {"x": x, "h": h}
        if case["grad"]:
            names = [k for k in ("x", "y", "weight", "post", "gate", "scale")
                     if isinstance(s[k], torch.Tensor)]
            grads = torch.autograd.grad((x, h), [s[k] for k in names], (s["d_x"], s["d_h"]))
            out |= {"d_" + k: g for k, g in zip(names, grads)}
        return out
    return {"update": ops.orthogonalize(s["g"], steps=_STEPS, coefficients=_QUINTIC, eps=_NS_EPS)}


@torch.no_grad()
def _run_plain(s):
    case = s["case"]
    dt = _DTYPES[case["dtype"]]
    if case["op"] == "logprobs":
        x = s["logits"].float()
        tokens = s["tokens"]
        live = tokens != _IGNORE
        d = x - x.amax(-1, keepdim=True)
        logz = d.exp().sum(-1, keepdim=True).log()
        lp = d - logz
        p = lp.exp()
        entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
        safe = torch.where(live, tokens, torch.zeros_like(tokens))[..., None]
        logp = torch.where(live, lp.gather(-1, safe)[..., 0], torch.zeros_like(entropy))
        out = {"logp": logp, "entropy": entropy}
        if case["top"]:
            order = x.sort(dim=-1, descending=True, stable=True).indices[..., :case["top"]]
            out |= {"top_logp": lp.gather(-1, order), "top_tokens": order.contiguous()}
        if case["grad"]:
            g = torch.where(live, s["d_logp"], torch.zeros_like(s["d_logp"]))[..., None]
            inner = torch.where(p > 0, lp, torch.zeros_like(lp)) + entropy[..., None]
            dx = -p * (g + s["d_entropy"][..., None] * inner)
            dx.scatter_add_(-1, safe, g)
            out["d_logits"] = dx.to(dt)
        return out
    if case["op"] == "embed":
        w, tokens = s["weight"], s["tokens"]
        out = {"h": (w[tokens].float() * s["scale"]).to(dt)}
        if case["grad"]:
            dw = torch.zeros(w.shape, device=w.device, dtype=torch.float32)
            dw.index_add_(0, tokens, s["d_out"].float() * s["scale"])
            if case["padding"]:
                dw[0] = 0
            out["d_weight"] = dw.to(dt)
        return out
    if case["op"] == "norm":
        D = case["width"]
        y = s["y"].float()
        one = torch.ones((), device=y.device)
        z, ry = y, None
        if case["post"]:
            ry = torch.rsqrt(y.square().mean(-1, keepdim=True) + _NORM_EPS)
            z = y * ry * s["post"]
        gate = torch.sigmoid(s["gate"].float()) if case["gate"] else one
        scale = one if s["scale"] is None else s["scale"]
        xn = (s["x"].float() + scale * gate * z).to(dt)
        t = xn.float()
        rx = torch.rsqrt(t.square().mean(-1, keepdim=True) + _NORM_EPS)
        out = {"x": xn, "h": (t * rx * s["weight"]).to(dt)}
        if case["grad"]:
            dh = s["d_h"].float()
            gw = dh * s["weight"]
            dt_ = s["d_x"].float() + rx * gw - t * (rx ** 3) * (gw * t).sum(-1, keepdim=True) / D
            dz = dt_ * scale * gate
            dy = dz
            if case["post"]:
                pw = dz * s["post"]
                dy = ry * pw - y * (ry ** 3) * (pw * y).sum(-1, keepdim=True) / D
            out |= {"d_x": dt_.to(dt), "d_y": dy.to(dt), "d_weight": (dh * t * rx).sum(0)}
            if case["post"]:
                out["d_post"] = (dz * y * ry).sum(0)
            if case["gate"]:
                out["d_gate"] = (dt_ * scale * z * gate * (1 - gate)).to(dt)
            if case["scale"] == "vector":
                out["d_scale"] = (dt_ * gate * z).sum(0)
        return out
    g = s["g"].float()
    tall = case["m"] > case["n"]
    x = g.mT if tall else g
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + _NS_EPS)
    a, b, c = _QUINTIC
    for _ in range(_STEPS):
        A = x @ x.mT
        x = a * x + (b * A + c * (A @ A)) @ x
    return {"update": (x.mT if tall else x).contiguous().to(torch.bfloat16)}


# ------------------------------------------------------- definitions, 64 bits
def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "logprobs":
        rows = case["batch"] * case["tokens"]
        n = rows * case["vocab"]
        nbytes = n * e + rows * (8 + 8 + 12 * case["top"])
        flops = 6 * n
        if case["grad"]:
            nbytes += n * e + rows * 8
            flops += 7 * n
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "embed":
        N, V, D = case["count"], case["vocab"], case["width"]
        # tokens, one table row in for each distinct id (at most one per token), one row out
        nbytes = 8 * N + min(N, V) * D * e + N * D * e
        flops = N * D
        if case["grad"]:
            nbytes += N * D * e + V * D * e
            flops += 2 * N * D
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "norm":
        n, D = case["rows"] * case["width"], case["width"]
        tensors = 4 + case["gate"]
        flops = 10 * n
        if case["grad"]:
            tensors += 4 + case["gate"]
            flops += 20 * n
        return {"bytes": tensors * n * e + 16 * D, "flops": flops}
    L, m, n = case["count"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # the two symmetric products need half their entries
    per = m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n
    return {"bytes": L * m * n * (e + 2), "flops": L * _STEPS * per}


@torch.no_grad()
def exact(case, seed):
    s = prepare(case, seed)
    f64 = torch.float64
    if case["op"] == "logprobs":
        B, T, V, k = case["batch"], case["tokens"], case["vocab"], case["top"]
        logits = s["logits"].detach()
        rows = {"logp": [], "entropy": [], "top_logp": [], "top_tokens": [], "d_logits": []}
        # blocks of positions keep the 64-bit temporaries small
        step = max(1, (1 << 26) // (B * V))
        for t0 in range(0, T, step):
            x = logits[:, t0:t0 + step].to(f64)
            tok = s["tokens"][:, t0:t0 + step]
            lse = torch.logsumexp(x, -1)
            lp = x - lse[..., None]
            p = lp.exp()
            plp = torch.nan_to_num(p * lp, nan=0.0)
            H = -plp.sum(-1)
            live = (tok != _IGNORE)
            hit = torch.zeros_like(x).scatter_(-1, tok.clamp(min=0)[..., None], 1.0)
            hit = hit * live[..., None].to(f64)
            picked = torch.nan_to_num(x, neginf=0.0) * hit
            rows["logp"].append(picked.sum(-1) - lse * live)
            rows["entropy"].append(H)
            if k:
                # one extreme at a time, the lowest index among equals
                left = x.clone()
                ids = []
                at = torch.arange(V, device=x.device)
                for _ in range(k):
                    best = left.amax(-1, keepdim=True)
                    i = torch.where(left == best, at, V).amin(-1, keepdim=True)
                    ids.append(i)
                    left.scatter_(-1, i, -math.inf)
                ids = torch.cat(ids, -1)
                rows["top_tokens"].append(ids)
                rows["top_logp"].append(lp.gather(-1, ids))
            if case["grad"]:
                g = s["d_logp"][:, t0:t0 + step].to(f64)[..., None]
                dH = s["d_entropy"][:, t0:t0 + step].to(f64)[..., None]
                rows["d_logits"].append(g * (hit - p * live[..., None]) - dH * (plp + p * H[..., None]))
        out = {}
        for name in ("logp", "entropy") + (("top_logp", "top_tokens") if k else ()) + \
                (("d_logits",) if case["grad"] else ()):
            out[name] = torch.cat(rows[name], 1)
        return out
    if case["op"] == "embed":
        w, tokens = s["weight"].detach(), s["tokens"]
        out = {"h": torch.index_select(w, 0, tokens).to(f64) * s["scale"]}
        if case["grad"]:
            dw = torch.zeros(w.shape, device=w.device, dtype=f64)
            live = tokens != 0 if case["padding"] else torch.ones_like(tokens, dtype=torch.bool)
            dw.index_put_((tokens[live],), s["d_out"][live].to(f64), accumulate=True)
            out["d_weight"] = dw * s["scale"]
        return out
    if case["op"] == "norm":
        # the residual stream is kept in its own type: that rounding is part of the operator
        y = s["y"].detach().to(f64)
        D = case["width"]
        full = {k: (v.detach().to(f64) if isinstance(v, torch.Tensor) else v) for k, v in s.items()}
        ny = (y.pow(2).sum(-1, keepdim=True) / D + _NORM_EPS).sqrt() if case["post"] else None
        yh = y / ny if case["post"] else y
        z = yh * full["post"] if case["post"] else yh
        sg = 1 / (1 + torch.exp(-full["gate"])) if case["gate"] else torch.ones_like(y)
        sc = 1.0 if full["scale"] is None else full["scale"]
        xs = full["x"] + sc * sg * z
        t = xs.to(torch.float32).to(_DTYPES[case["dtype"]]).to(f64)
        nt = (t.pow(2).sum(-1, keepdim=True) / D + _NORM_EPS).sqrt()
        th = t / nt
        out = {"x": xs, "h": th * full["weight"]}
        if case["grad"]:
            dth = full["d_h"] * full["weight"]
            dt = full["d_x"] + (dth - th * (dth * th).sum(-1, keepdim=True) / D) / nt
            dz = dt * (sc * sg)
            if case["post"]:
                dyh = dz * full["post"]
                dy = (dyh - yh * (dyh * yh).sum(-1, keepdim=True) / D) / ny
            else:
                dy = dz
            out |= {"d_x": dt, "d_y": dy, "d_weight": torch.einsum("nd,nd->d", full["d_h"], th)}
            if case["post"]:
                out["d_post"] = torch.einsum("nd,nd->d", dz, yh)
            if case["gate"]:
                out["d_gate"] = dt * sc * z * (sg - sg * sg)
            if case["scale"] == "vector":
                out["d_scale"] = torch.einsum("nd,nd->d", dt, sg * z)
        return out
    g = s["g"].to(f64)
    x = g / (torch.linalg.matrix_norm(g)[..., None, None] + _NS_EPS)
    a, b, c = _QUINTIC
    eye = torch.eye(min(case["m"], case["n"]), device=g.device, dtype=f64)
    for _ in range(_STEPS):
        # the polynomial of the smaller Gram matrix, from whichever side that is
        if case["m"] > case["n"]:
            G = x.mT @ x
            x = torch.matmul(x, a * eye + torch.matmul(G, b * eye + c * G))
        else:
            G = x @ x.mT
            x = torch.matmul(a * eye + torch.matmul(G, b * eye + c * G), x)
    return {"update": x}

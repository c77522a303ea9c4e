"""The language-model operators in the paths that call them: a training step of the
model with the embedding, residual norms and loss as libcyfa operators and Muon as
the optimizer, scoring, and the graph decoder's ratings."""

import math

import pytest
import torch

from gpu_util import rel_l2, seeded
from oracle import cyfa_oracle as O

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)


def _model(seed=0):
    from cyclic_flow_attention.models.cyfa import CyclicFlowAttentionConfig
    from cyclic_flow_attention.utils import initialize_model

    cfg = CyclicFlowAttentionConfig(hidden_size=256, num_heads=2, head_dim=128,
                                    num_hidden_layers=2, vocab_size=512)
    m = initialize_model(cfg, generator=seeded(seed))
    with torch.no_grad():
        for blk in m.model.layers:
            blk.attn.readout.add_(0.05 * torch.randn(blk.attn.readout.shape, generator=seeded(1)))
    return cfg, m.cuda().train()


def _grads(m, ids, labels):
    m.zero_grad(set_to_none=True)
    out = m(ids, labels=labels)
    out["loss"].backward()
    return out["loss"].detach(), {n: p.grad.detach().clone() for n, p in m.named_parameters()}


def test_fused_step_matches_the_glue_step():
    """Same weights and batch: the loss of both paths is the same fp32 sum in another
    order (2^-20 relative), and each gradient of the fused path is no further from
    the fp32 oracle's than the PyTorch glue's, up to the rounding of one bf16 step.
    Both are the same bf16 computation with roundings in other places, so their
    errors are two draws of one noise: its norm is compared where it averages over
    1000 entries or more (to a few percent), and over all parameters together; the
    gate parameters' gradients, a few cancelling sums each, say nothing alone."""
    cfg, m = _model()
    ids = torch.randint(0, cfg.vocab_size, (2, 160), generator=seeded(3)).cuda()
    labels = ids.clone()
    labels[0, 100:] = -100
    loss0, g0 = _grads(m, ids, labels)
    loss1, g1 = _grads(m.fuse_training(), ids, labels)
    loss2, g2 = _grads(m.fuse_training(False), ids, labels)
    assert torch.equal(loss0, loss2) and all(torch.equal(g0[n], g2[n]) for n in g0)
    params = {n: t.detach().float().cpu().requires_grad_() for n, t in m.named_parameters()}
    logits = O.cyfa_lm(params, ids.cpu(), cfg.num_hidden_layers, cfg.num_heads, cfg.head_dim,
                       cfg.head_dim)
    ref = torch.nn.functional.cross_entropy(logits[:, :-1].reshape(-1, cfg.vocab_size),
                                            labels[:, 1:].reshape(-1).cpu(), ignore_index=-100)
    ref.backward()
    # both paths make the same bf16 logits up to single roundings
    assert abs(float(loss1) - float(loss0)) < 2.0 ** -8 * abs(float(loss0))
    for n, p in params.items():
        e0, e1 = rel_l2(g0[n], p.grad), rel_l2(g1[n], p.grad)
        assert g1[n].dtype == g0[n].dtype
        assert p.numel() < 1000 or e1 < 1.2 * e0 + 2.0 ** -8, (n, e0, e1)
    whole = [torch.cat([d[n].float().cpu().reshape(-1) for n in params]) for d in (g0, g1)]
    ref = torch.cat([p.grad.reshape(-1) for p in params.values()])
    assert rel_l2(whole[1], ref) < 1.2 * rel_l2(whole[0], ref)


def test_fused_step_with_a_padded_batch():
    """A right-padded batch with its attention mask, and one row without any label:
    both paths are one bf16 computation rounded in other places, at most 40 roundings
    of 2^-8 one after the other between a parameter's gradient and the inputs."""
    cfg, m = _model(4)
    ids = torch.randint(0, cfg.vocab_size, (3, 130), generator=seeded(5)).cuda()
    mask = torch.ones_like(ids)
    mask[0, 77:] = 0
    labels = ids.masked_fill(mask == 0, -100)
    labels[2] = -100
    got = []
    for on in (False, True):
        m.fuse_training(on).zero_grad(set_to_none=True)
        loss = m(ids, labels=labels, attention_mask=mask)["loss"]
        loss.backward()
        got.append((loss.detach(), torch.cat([p.grad.float().reshape(-1) for p in m.parameters()])))
    assert abs(float(got[1][0]) - float(got[0][0])) < 2.0 ** -8 * abs(float(got[0][0]))
    assert rel_l2(got[1][1], got[0][1]) < 40 * 2.0 ** -8


def test_fused_step_captured_and_repeated():
    """The fused forward and backward in one CUDA graph, replayed: the same gradients
    as eager, bit for bit (no atomics anywhere)."""
    from cyclic_flow_attention.graphs import GraphedStep

    cfg, m = _model()
    m.fuse_training()
    ids = torch.randint(0, cfg.vocab_size, (2, 128), generator=seeded(4)).cuda()
    loss, g = _grads(m, ids, ids)
    again, h = _grads(m, ids, ids)
    assert torch.equal(loss, again) and all(torch.equal(g[n], h[n]) for n in g)
    del loss, again, h
    params = [p for p in m.parameters()]

    def step(x):
        out = m(x, labels=x)["loss"]
        out.backward()
        return out.detach()

    captured = GraphedStep(step, [ids.clone()], params=params)
    other = torch.randint(0, cfg.vocab_size, (2, 128), generator=seeded(5)).cuda()
    captured(other)
    captured(ids)
    for (n, p) in m.named_parameters():
        assert torch.equal(p.grad, g[n]), n


def test_score_matches_log_softmax():
    cfg, m = _model()
    m.eval()
    ids = torch.randint(0, cfg.vocab_size, (3, 96), generator=seeded(6)).cuda()
    mask = torch.ones_like(ids)
    mask[1, 70:] = 0
    r = m.score(ids, mask, top=4)
    with torch.no_grad():
        hidden, _ = m.model(ids, None, False, mask)
        lp = torch.log_softmax(m.lm_head(hidden)[:, :-1].double(), -1)
    want = lp.gather(-1, ids[:, 1:, None])[..., 0]
    live = mask[:, 1:] == 1
    assert (r.logp.double() - want)[live].abs().max() < 2.0 ** -15
    assert (r.logp[~live] == 0).all()
    assert (r.entropy.double() + (lp.exp() * lp).sum(-1))[live].abs().max() < 2.0 ** -14
    assert torch.equal(r.top_tokens[live], lp.sort(dim=-1, descending=True, stable=True)
                       .indices[..., :4][live])


def test_graphed_decoder_scores():
    from cyclic_flow_attention.generation import GraphedDecoder

    cfg, m = _model()
    m.eval()
    ids = torch.randint(0, cfg.vocab_size, (4, 64), generator=seeded(7)).cuda()
    plain = GraphedDecoder(m).generate(ids, 6)
    dec = GraphedDecoder(m, top=3)
    tokens = [dec.prefill(ids)]
    with torch.no_grad():
        logits, cache = m.model(ids, use_cache=True)
        logits = m.lm_head(logits[:, -1])
        for step in range(6):
            if step:
                tokens.append(dec.step().clone())
                logits, cache = m.decode_step(tokens[step - 1], cache)
            s = dec.scores
            lp = torch.log_softmax(logits.double(), -1)
            assert (s.logp.double() - lp.gather(-1, tokens[step])[:, 0]).abs().max() < 2.0 ** -15
            assert torch.equal(s.top_tokens[:, :1], tokens[step])
            assert torch.equal(s.top_tokens, lp.sort(dim=-1, descending=True, stable=True)
                               .indices[:, :3])
    assert torch.equal(torch.cat(tokens, 1), plain)
    assert GraphedDecoder(m).scores is None


def _ns(g, steps=5):
    x = g.double()
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    x = x / (x.norm() + 1e-7)
    for _ in range(steps):
        A = x @ x.T
        x = QUINTIC[0] * x + (QUINTIC[1] * A + QUINTIC[2] * A @ A) @ x
    return x.T if tall else x


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_matches_the_formula(nesterov):
    """Three steps of mixed parameters against 64 bits.  A step's update is off by its
    rounding to bf16 (2^-8 relative) times lr; masters by fp32 roundings besides."""
    from training.optim import AdamW, Muon

    torch.manual_seed(0)
    shapes = [("a.weight", (96, 200)), ("b.weight", (200, 96)), ("c.weight", (96, 200)), ("d.bias", (33,)),
              ("embeddings.weight", (50, 40)), ("e.weight", (5, 7)), ("r", (2, 9, 9))]
    dts = [torch.bfloat16, torch.float32, torch.bfloat16, torch.float32, torch.bfloat16, torch.float32,
           torch.float32]
    ps = [(n, torch.randn(s, device="cuda").to(dt).requires_grad_()) for (n, s), dt in zip(shapes, dts)]
    lr, mu, wd = 0.02, 0.9, 0.1
    opt = Muon(ps, lr=lr, momentum=mu, nesterov=nesterov, weight_decay=wd, adamw_lr=1e-3)
    ref_ps = [(n, p.detach().clone().requires_grad_()) for n, p in ps]
    others = AdamW([q for q in ref_ps if q[1].dim() != 2 or "embeddings" in q[0]], lr=1e-3)
    master = {n: p.detach().double() for n, p in ps}
    mom = {n: torch.zeros_like(w) for n, w in master.items()}
    assert [g.get("matrix", False) for g in opt.param_groups] == [True, False]
    for step in range(3):
        gs = [torch.randn(p.shape, device="cuda").to(p.dtype) for _, p in ps]
        for (_, p), (_, q), g in zip(ps, ref_ps, gs):
            p.grad, q.grad = g, g.clone()
        opt.accumulate_param_grads()
        others.accumulate_param_grads()
        opt.step()
        others.step()
        for (n, p), g in zip(ps, gs):
            if p.dim() == 2 and "embeddings" not in n:
                mom[n] = mu * mom[n] + g.double()
                u = g.double() + mu * mom[n] if nesterov else mom[n]
                o = _ns(u)
                f = lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1]))
                master[n] = master[n] * (1 - lr * wd) - f * o
                got = {k: w for gr in opt.param_groups for k, w in zip(gr["names"], gr["master"])}[n]
                err = (got.double() - master[n]).norm() / (f * o.norm() * (step + 1))
                assert err < 2.0 ** -8, (n, step, float(err))
                assert torch.equal(p.detach(), got.to(p.dtype))
                master[n] = got.double()
    for (n, p), (_, q) in zip(ps, ref_ps):
        if p.dim() != 2 or "embeddings" in n:
            assert torch.equal(p.detach(), q.detach()), n


def test_whole_training_step():
    """Embedding, residual norms, loss and Muon together, as a program uses them: three
    steps with clipping leave every parameter finite and changed."""
    from training.optim import Muon

    cfg, m = _model()
    m.fuse_training()
    before = {n: p.detach().clone() for n, p in m.named_parameters()}
    opt = Muon(m.named_parameters(), lr=0.01)
    matrices = opt.param_groups[0]["names"]
    assert any("down_proj" in n for n in matrices) and not any("embeddings" in n for n in matrices)
    ids = torch.randint(0, cfg.vocab_size, (2, 128), generator=seeded(8)).cuda()
    for _ in range(3):
        opt.backward(m(ids, labels=ids)["loss"])
        assert torch.isfinite(opt.clip_grad_norm(1.0))
        opt.step()
    for n, p in m.named_parameters():
        assert torch.isfinite(p).all() and not torch.equal(p.detach(), before[n]), n


def test_second_derivatives_are_refused():
    """A gradient taken with create_graph has the ordinary values; differentiating it
    again is an error, not a silent zero."""
    from cyclic_flow_attention.ops import embed_tokens, residual_norm, token_log_probs

    x = torch.randn(6, 32, device="cuda", requires_grad=True)
    w = torch.rand(32, device="cuda", requires_grad=True)
    t = torch.tensor([3, 1, 3, 0, 5, 5], device="cuda")
    for f, saved in ((lambda: residual_norm(x, x, w)[1], True),
                     (lambda: token_log_probs(x, t).logp, True), (lambda: embed_tokens(t, x), False)):
        d = torch.randn_like(f())
        plain, = torch.autograd.grad(f(), x, d)
        for given in (d, d.clone().requires_grad_()):
            g, = torch.autograd.grad(f(), x, given, create_graph=True)
            assert torch.equal(g, plain)
            for source, on in ((x, saved), (given, given.requires_grad)):
                if on:
                    with pytest.raises(RuntimeError, match="second derivative"):
                        torch.autograd.grad(g.sum(), source, retain_graph=True)
